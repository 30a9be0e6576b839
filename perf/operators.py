"""Performance cases of a speculative decoding step on the packed KV cache: several drafted tokens of a sequence, arranged
as a tree, go through the model at once, are attended against the cache, verified, and the accepted ones stay.

A case is a dict of plain values; `kind` picks the call:

  write    ops.KVCache.write_qkv (QKV projection -> normed, rotated queries; keys and values into the cache)
  attend   ops.KVCache.attend_tree (the nodes of a tree against the cache and their own ancestors)
  verify   ops.verify_tree (which drafted tokens stay, and the token behind them)
  keep     ops.KVCache.keep (the accepted nodes' rows move together)

`own` chooses between these calls and their plain forms in elementary torch operations.  `exact` has the computed results
in 64 bits, from the raw inputs, with its own quantiser and rotation.  Inputs are synthetic: activations, keys and values
~ N(0, 1) in bf16, a few key channels larger than the rest; distributions over the vocabulary are softmaxes of normal
logits, the drafts' those of the same logits with noise.
"""

import math

import torch

from ms_kernel_b200 import ops

own = False

DEV = "cuda"
GS = 2                      # the group size of every configuration of this repository
D = 128                     # head dimension of every configuration of this repository
NB = D // 32
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a short conversation, a small tree: the smallest attention call, launch latency counts
        {"name": "attend 32/8 B1 T8 509", "kind": "attend", "B": 1, "T": 8, "Hq": 32, "Hkv": 8, "ctx": 509, "u": 4},
        # one long conversation with a large odd tree, eight query heads to a key head
        {"name": "attend 64/8 B1 T61 16381", "kind": "attend", "B": 1, "T": 61, "Hq": 64, "Hkv": 8, "ctx": 16381, "u": 4},
        # many long conversations of different lengths: the largest attention call
        {"name": "attend 32/8 B16 T16 32752", "kind": "attend", "B": 16, "T": 16, "Hq": 32, "Hkv": 8, "ctx": 32752, "u": 4},
        # three query heads to a key head, the 5+3 bit format, a handful of sequences
        {"name": "attend 24/8 B5 T7 4099 u3", "kind": "attend", "B": 5, "T": 7, "Hq": 24, "Hkv": 8, "ctx": 4099, "u": 3},
        # ordinary decoding of one token: the smallest write
        {"name": "write 32/8 B1 T1", "kind": "write", "B": 1, "T": 1, "Hq": 32, "Hkv": 8, "Lcap": 4096, "u": 4, "tree": False},
        # the prompt of one conversation, of odd length
        {"name": "write 32/8 B1 T8191", "kind": "write", "B": 1, "T": 8191, "Hq": 32, "Hkv": 8, "Lcap": 8192, "u": 4, "tree": False},
        # drafted trees of a batch: positions by depth, sequences at different slots, some trees smaller than others
        {"name": "write 32/8 B16 T16 tree", "kind": "write", "B": 16, "T": 16, "Hq": 32, "Hkv": 8, "Lcap": 2048, "u": 4, "tree": True},
        # one sequence, drafts taken as they are (no draft distribution)
        {"name": "verify B1 T8 V32000", "kind": "verify", "B": 1, "T": 8, "V": 32000, "drafts": False},
        # a batch with large trees drawn from a draft model's distributions
        {"name": "verify B16 T64 V128256", "kind": "verify", "B": 16, "T": 64, "V": 128256, "drafts": True},
        # the accepted nodes of one small tree
        {"name": "keep B1 T8", "kind": "keep", "B": 1, "T": 8, "Hkv": 8, "Lcap": 1024, "u": 4},
        # the same after a batch with large trees
        {"name": "keep B64 T61", "kind": "keep", "B": 64, "T": 61, "Hkv": 8, "Lcap": 1024, "u": 4},
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """Trees of 2 to 64 nodes over contexts of 16 to 32752 keys, one to eight query heads to a key head, batches of 1 to 16
    (64 where only the cache is touched), any u; writes of one token to a prompt of 8191; vocabularies of 1000 to 128256."""
    kind = rng.choice(["attend"] * 4 + ["write"] * 3 + ["verify"] * 2 + ["keep"])
    u = rng.choice([4, 4, 3, 2])
    if kind == "attend":
        Hkv, G, T = rng.choice([1, 2, 4, 8]), rng.randint(1, 8), _log_int(rng, 2, 64)
        B = _log_int(rng, 1, 16)
        most = 16 * 8 * 32752 * 64 // (B * Hkv * max(64, T * G))
        return {"kind": kind, "B": B, "T": T, "Hq": Hkv * G, "Hkv": Hkv, "ctx": _log_int(rng, 16, min(32752, most)), "u": u}
    if kind == "write":
        Hkv, G, tree = rng.choice([1, 2, 4, 8]), rng.randint(1, 8), rng.random() < 0.5
        B = _log_int(rng, 1, 16)
        T = _log_int(rng, 2, 64) if tree else rng.choice([1, _log_int(rng, 2, 8191 // B)])
        return {"kind": kind, "B": B, "T": T, "Hq": Hkv * G, "Hkv": Hkv, "Lcap": _log_int(rng, T + 1, max(2048, T + 65)), "u": u, "tree": tree}
    if kind == "verify":
        return {"kind": kind, "B": _log_int(rng, 1, 16), "T": _log_int(rng, 2, 64), "V": _log_int(rng, 1000, 128256),
                "drafts": rng.random() < 0.6}
    return {"kind": kind, "B": _log_int(rng, 1, 64), "T": _log_int(rng, 2, 64), "Hkv": rng.choice([1, 2, 4, 8]),
            "Lcap": _log_int(rng, 128, 1024), "u": u}


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 64 + stream)


def _cpu_gen(seed, stream):
    return torch.Generator().manual_seed(int(seed) * 64 + stream)


def _randn(shape, gen):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.bfloat16)


def _keys_values(B, Hkv, L, seed):
    g = _gen(seed, 1)
    K, V = _randn((B, Hkv, L, D), g), _randn((B, Hkv, L, D), g)
    K[..., 5] *= 4                                       # keys have a few channels that are larger than the rest
    K[..., 77] *= 3
    return K, V


def _parents(B, T, seed):
    """Random trees: every node hangs on the one before it or on any earlier one."""
    g = _cpu_gen(seed, 2)
    any_of = (torch.rand((B, T), generator=g) * torch.arange(T).clamp_min(1)).long()
    before = torch.arange(T).expand(B, T) - 1
    par = torch.where(torch.rand((B, T), generator=g) < 0.5, before, any_of)
    par[:, 0] = -1
    return par.to(torch.int32)


def _masks_depths(parents):
    """Bit j of mask[b, i]: node i sees node j (itself and its ancestors); depth below the root."""
    B, T = parents.shape
    par = parents.tolist()
    mask, depth = [[0] * T for _ in range(B)], [[0] * T for _ in range(B)]
    for b in range(B):
        for i in range(T):
            p = par[b][i]
            mask[b][i] = (1 << i) | (mask[b][p] if p >= 0 else 0)
            depth[b][i] = depth[b][p] + 1 if p >= 0 else 0
    signed = [[m - (1 << 64) if m >> 63 else m for m in row] for row in mask]
    return torch.tensor(signed, dtype=torch.int64), torch.tensor(depth, dtype=torch.int32)


def _lens(B, most, seed):
    """Ragged lengths of a batch (the longest is `most`)."""
    f = torch.rand(B, generator=_cpu_gen(seed, 3))
    lens = (most * (0.5 + 0.5 * f)).to(torch.int32).clamp(0, most)
    lens[0] = most
    return lens


def _rope_tables(rows):
    inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device=DEV).double() / D))
    f = torch.outer(torch.arange(rows, device=DEV).double(), inv)
    return torch.cos(f).float().contiguous(), torch.sin(f).float().contiguous()


def _capacity(L):
    return (L + 15) // 16 * 16


def _attend_inputs(case, seed):
    B, T = case["B"], case["T"]
    q = _randn((B, T, case["Hq"], D), _gen(seed, 4))
    mask, _ = _masks_depths(_parents(B, T, seed))
    return q, mask.to(DEV), _lens(B, case["ctx"], seed)


def _write_inputs(case, seed):
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    g = _gen(seed, 5)
    qkv = _randn((B, T, (Hq + 2 * Hkv) * D), g)
    gains = [(1.0 + 0.25 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2)]
    start = _lens(B, case["Lcap"] - T, seed)
    pos = counts = None
    if case["tree"]:
        _, depth = _masks_depths(_parents(B, T, seed))
        pos = (start[:, None] + depth).to(torch.int32).to(DEV)
        counts = _lens(B, T, seed + 1).clamp_min(1).to(DEV)
    return qkv, gains[0], gains[1], start.to(DEV), pos, counts


def _verify_inputs(case, seed):
    B, T, V = case["B"], case["T"], case["V"]
    g = _gen(seed, 6)
    target = torch.empty((B, T, V), device=DEV)
    draft = torch.empty((B, T, V), device=DEV) if case["drafts"] else None
    likely = torch.empty((B, T, T), dtype=torch.int64, device=DEV)
    for b in range(B):
        z = 3.0 * torch.randn((T, V), generator=g, device=DEV)
        target[b] = torch.softmax(z, -1)
        z += 0.7 * torch.randn((T, V), generator=g, device=DEV)
        z = torch.softmax(z, -1)
        if case["drafts"]:
            draft[b] = z
            likely[b] = torch.multinomial(z, T, replacement=True, generator=g)
        else:
            likely[b] = torch.topk(z, T).indices
    parents = _parents(B, T, seed).to(DEV)
    # a node's token comes from its parent's row; siblings take different columns of `likely`
    row = likely.gather(1, parents.long().clamp_min(0)[..., None].expand(B, T, T))
    same = (parents[:, :, None] == parents[:, None, :]) & torch.ones((T, T), dtype=torch.bool, device=DEV).tril(-1)
    tokens = row.gather(2, same.sum(-1)[..., None])[..., 0].to(torch.int32)
    return target, draft, tokens, parents, torch.rand((B, T), generator=g, device=DEV)


def _keep_inputs(case, seed):
    """For each sequence a way down a tree: ascending node numbers that begin with the root."""
    B, T = case["B"], case["T"]
    par = _parents(B, T, seed).tolist()
    pick = torch.randint(0, T, (B,), generator=_cpu_gen(seed, 7)).tolist()
    path, count = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        way, i = [], pick[b]
        while i >= 0:
            way.append(i)
            i = par[b][i]
        way.reverse()
        path[b, : len(way)] = torch.tensor(way, dtype=torch.int32)
        count[b] = len(way)
    return _lens(B, case["Lcap"] - T, seed).to(DEV), path.to(DEV), count.to(DEV)


def prepare(case, seed):
    kind = case["kind"]
    if kind == "verify":
        target, draft, tokens, parents, uniforms = _verify_inputs(case, seed)
        return {"kind": kind, "target": target, "draft": draft, "tokens": tokens, "parents": parents, "uniforms": uniforms}
    B, T, Hkv, u = case["B"], case["T"], case["Hkv"], case["u"]
    if kind == "attend":
        Lk = case["ctx"] + T
        cache = ops.KVCache(B, Hkv, D, _capacity(Lk), u, GS, DEV)
        cache.fill(*_keys_values(B, Hkv, Lk, seed))
        q, mask, lens = _attend_inputs(case, seed)
        return {"kind": kind, "cache": cache, "q": q, "mask": mask, "lens": lens.to(DEV), "Lk": Lk}
    cache = ops.KVCache(B, Hkv, D, case["Lcap"], u, GS, DEV)
    if kind == "write":
        qkv, qg, kg, start, pos, counts = _write_inputs(case, seed)
        return {"kind": kind, "cache": cache, "Hq": case["Hq"], "qkv": qkv, "q_gain": qg, "k_gain": kg, "start": start, "pos": pos,
                "counts": counts, "rope": _rope_tables(case["Lcap"])}
    cache.fill(*_keys_values(B, Hkv, case["Lcap"], seed))
    start, path, count = _keep_inputs(case, seed)
    return {"kind": kind, "cache": cache, "start": start, "path": path, "count": count}


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["kind"]
    if kind == "verify":
        if own:
            return list(ops.verify_tree(state["target"], state["tokens"], state["parents"], state["uniforms"], state["draft"]))
        return _plain_verify(state)
    c = state["cache"]
    if kind == "attend":
        if own:
            return c.attend_tree(state["q"], state["mask"], state["Lk"], state["lens"])
        return _plain_attend(state)
    if kind == "write":
        if own:
            q = c.write_qkv(state["qkv"], state["Hq"], state["start"], state["rope"], state["q_gain"], state["k_gain"], EPS,
                            pos=state["pos"], counts=state["counts"])
        else:
            q = _plain_write(state)
        return [q, *c.k, *c.v]
    if own:
        c.keep(state["start"], state["path"], state["count"])
    else:
        _plain_keep(state)
    return [*c.k, *c.v]


# ---------------------------------------------------------------------------------------------- plain forms
def _fields(plane, width, count):
    """Bytes [..., n] of a dense little-endian run of `count` two's-complement fields -> int16 [..., count]."""
    bits = (plane[..., None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1
    bits = bits.reshape(*plane.shape[:-1], -1)[..., : count * width].reshape(*plane.shape[:-1], count, width)
    weight = [1 << k for k in range(width)]
    weight[-1] = -weight[-1]
    return (bits.to(torch.float16) * torch.tensor(weight, device=DEV, dtype=torch.float16)).sum(-1)


def _run_of(codes, width):
    """Whole numbers [..., count] -> bytes of the dense little-endian run of their low `width` bits."""
    bits = (codes[..., None].to(torch.int32) >> torch.arange(width, device=DEV, dtype=torch.int32)) & 1
    bits = bits.reshape(*codes.shape[:-1], -1, 8)
    return (bits * (1 << torch.arange(8, device=DEV, dtype=torch.int32))).sum(-1).to(torch.uint8)


def _dequantised(planes, u):
    """Planes of one cache -> its values [B, Hkv, Lcap, D] in 32 bits."""
    e, upper, shared = planes
    up, sh = _fields(upper, 8 - u, 32), _fields(shared, u, 32 // GS)
    q = (up * (1 << u) + sh.repeat_interleave(GS, -1)).float()
    x = q * torch.exp2(e.float())[..., None]
    return x.permute(0, 1, 3, 2, 4).reshape(e.shape[0], e.shape[1], e.shape[3], D)


def _rotated(x):
    """The orthonormal Hadamard rotation of the last axis in 32 bits, stage by stage."""
    y, h = x.float(), 1
    while h < D:
        z = y.reshape(*x.shape[:-1], D // (2 * h), 2, h)
        y = torch.stack((z[..., 0, :] + z[..., 1, :], z[..., 0, :] - z[..., 1, :]), -2).reshape(x.shape)
        h *= 2
    return y * torch.tensor(1.0 / math.sqrt(D), dtype=torch.float32, device=DEV)


def _plain_attend(state):
    c, q, mask, lens = state["cache"], state["q"], state["mask"], state["lens"]
    B, T, Hq, _ = q.shape
    K, V = _dequantised(c.k, c.u), _dequantised(c.v, c.u)
    key = torch.arange(c.Lcap, device=DEV)
    node = key - lens[:, None]                                                       # [B, Lcap]
    bit = (mask[:, :, None] >> node.clamp(0, 63)[:, None]) & 1                       # [B, T, Lcap]
    seen = torch.where((node < 0)[:, None], True, (node < T)[:, None] & (bit == 1))
    G = Hq // c.Hkv
    qr = _rotated(q).reshape(B, T, c.Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, c.Hkv, T * G, D)
    s = torch.matmul(qr, K.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    s = s.reshape(B, c.Hkv, T, G, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).reshape(B, c.Hkv, T * G, -1)
    o = torch.matmul(p, V).reshape(B, c.Hkv, T, G, D).permute(0, 2, 1, 3, 4)
    return o.reshape(B, T, Hq, D).to(torch.bfloat16)


def _quantised(x, u):
    """x [..., D] -> exponent, upper and shared bytes of its 32-blocks: grid 2^(floor(log2 max|x|) - 6), upper codes on 2^u
    times the grid, one shared code for the mean residual of each pair; in 64 bits, where a value may lie on a half."""
    b = x.double().reshape(*x.shape[:-1], NB, 32)
    e = (torch.frexp(b.abs().amax(-1, keepdim=True).clamp_min(1e-30)).exponent - 7).clamp(-127, 127)
    fine = torch.exp2(e.double())
    up = torch.round(b / (fine * (1 << u))).clamp(-((1 << (7 - u)) - 1), (1 << (7 - u)) - 1)
    res = (b - up * fine * (1 << u)).reshape(*b.shape[:-1], 32 // GS, GS)
    sh = torch.round(res.sum(-1) / GS / fine).clamp(-(1 << (u - 1)), (1 << (u - 1)) - 1)
    return e[..., 0].to(torch.int8), _run_of(up, 8 - u), _run_of(sh, u)


def _normed(x, gain):
    """x [..., D] times the reciprocal root of its mean square, times gain; the mean in 64 bits, where the codes that follow
    may lie on a half."""
    x64 = x.double()
    r = torch.rsqrt(x64.square().mean(-1, keepdim=True) + EPS).float()
    return x.float() * r * gain.float()


def _plain_write(state):
    c, Hq, start, pos, counts = state["cache"], state["Hq"], state["start"], state["pos"], state["counts"]
    qkv = state["qkv"]
    B, T, _ = qkv.shape
    heads = qkv.reshape(B, T, Hq + 2 * c.Hkv, D)
    slot = start[:, None].long() + torch.arange(T, device=DEV)                       # [B, T]
    at = slot if pos is None else pos.long()
    y = torch.cat((_normed(heads[:, :, :Hq], state["q_gain"]), _normed(heads[:, :, Hq:Hq + c.Hkv], state["k_gain"])), 2)
    cos, sin = (t[at][:, :, None] for t in state["rope"])
    a, b = y[..., 0::2], y[..., 1::2]
    y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(y.shape).to(torch.bfloat16)
    live = torch.arange(T, device=DEV) < (T if counts is None else counts[:, None])
    live = live.expand(B, T)
    # in the place of padding the first token is written once more
    seq, dest = torch.arange(B, device=DEV)[:, None].expand(B, T), torch.where(live, slot, slot[:, :1])
    take = torch.where(live, torch.arange(T, device=DEV), 0)
    for X, planes in ((_rotated(y[:, :, Hq:]), c.k), (heads[:, :, Hq + c.Hkv:], c.v)):
        for code, plane in zip(_quantised(X, c.u), planes):                          # code [B, T, Hkv, NB, ...]
            plane.transpose(1, 3).transpose(2, 3)[seq, dest] = code[seq, take]
    return torch.where(live[:, :, None, None], y[:, :, :Hq], 0.0).to(torch.bfloat16)


def _positive(p):
    """Probabilities in 64 bits; what is not positive and finite counts as nothing."""
    p = p.double()
    return torch.where((p > 0) & (p < math.inf), p, 0.0)


def _plain_verify(state):
    target, draft, tokens, parents, u = (state[k] for k in ("target", "draft", "tokens", "parents", "uniforms"))
    B, T, V = target.shape
    rows = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.int64, device=DEV)
    path = torch.full((B, T), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    count = torch.ones(B, dtype=torch.int32, device=DEV)
    r, Z = _positive(target[:, 0]), torch.ones(B, dtype=torch.float64, device=DEV)
    place = torch.arange(T, device=DEV)
    for j in range(1, T):                                # the way down the tree depends on every decision before it
        x = tokens[:, j].long()
        child = (parents[:, j] == cur) & (x >= 0) & (x < V)
        x = x.clamp(0, V - 1)
        rx = r[rows, x]
        q = None if draft is None else _positive(draft[rows, cur])
        qx = 1.0 if draft is None else q[rows, x]
        accept = child & (u[:, j].double() * qx * Z < rx)
        reject = child & ~accept
        if draft is None:
            r[rows, x] = torch.where(reject, 0.0, rx)
            Z = torch.where(reject, Z - rx, Z)
        else:
            r = torch.where(reject[:, None], (r - Z[:, None] * q).clamp_min(0.0), r)
            Z = torch.where(reject, r.sum(-1), Z)
        path = torch.where(accept[:, None] & (place == count[:, None]), j, path)
        count = count + accept.to(torch.int32)
        cur = torch.where(accept, j, cur)
        r = torch.where(accept[:, None], _positive(target[:, j]), r)
        Z = torch.where(accept, 1.0, Z)
    r = torch.where((r.sum(-1) > 0)[:, None], r, _positive(target[rows, cur]))
    total = r.sum(-1)
    token = (r.cumsum(-1) <= (u[:, 0].double() * total)[:, None]).sum(-1)
    last = torch.where(r > 0, torch.arange(V, device=DEV), -1).amax(-1)
    return [path, count, torch.minimum(token, last).to(torch.int32)]


def _plain_keep(state):
    c, start, path, count = state["cache"], state["start"], state["path"], state["count"]
    B, T = path.shape
    k = torch.arange(T, device=DEV)
    stays = k < count[:, None]
    seq = torch.arange(B, device=DEV)[:, None].expand(B, T)
    dest = start[:, None].long() + k
    source = torch.where(stays, start[:, None].long() + path, dest)
    for plane in (*c.k, *c.v):
        by_slot = plane.transpose(1, 3).transpose(2, 3)                              # [B, Lcap, Hkv, NB, ...]
        by_slot[seq, dest] = by_slot[seq, source]


# ---------------------------------------------------------------------------------------------- what a pass needs
def _row_bytes(u):
    return NB * (32 * (8 - u) // 8 + 32 // GS * u // 8 + 1)                          # one packed row of a key or value head


def work(case):
    kind, B, T = case["kind"], case["B"], case["T"]
    if kind == "verify":
        b = B * case["V"] * 4 * (2 if case["drafts"] else 1) + 20 * B * T            # the last row visited, p and q
        return {"bytes": float(b), "flops": float(B * case["V"] * (3 if case["drafts"] else 1))}
    Hkv, row = case["Hkv"], _row_bytes(case["u"])
    if kind == "attend":
        keys = case["ctx"] * (0.75 * (B - 1) + 1) + B * T                            # of the whole batch
        return {"bytes": float(keys * Hkv * 2 * row + 4 * B * T * case["Hq"] * D), "flops": float(4 * keys * T * case["Hq"] * D)}
    if kind == "write":
        n = (0.75 * (B - 1) + 1) * T if case["tree"] else B * T
        heads = case["Hq"] + 2 * Hkv
        return {"bytes": float(n * (2 * D * (heads + case["Hq"]) + 2 * Hkv * row + 4 * D)), "flops": float(n * heads * D * 12)}
    return {"bytes": float(B * (T ** 0.5) * Hkv * 4 * row), "flops": 0.0}


# ---------------------------------------------------------------------------------------------- 64-bit results
def _hadamard64():
    """Sylvester's matrix of order D, orthonormal."""
    h = torch.ones((1, 1), dtype=torch.float64, device=DEV)
    while h.shape[0] < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / math.sqrt(D)


def _stored64(x, u):
    """The values that the cache stands for after x [L, D] was written to it."""
    b = x.double().reshape(-1, NB, 32)
    grid = torch.exp2((torch.frexp(b.abs().amax(-1, keepdim=True).clamp_min(1e-30)).exponent - 7).clamp(-127, 127).double())
    top = 2 ** (7 - u) - 1
    coarse = torch.round(b / grid / 2 ** u).clamp(-top, top) * 2 ** u
    left = (b / grid - coarse).reshape(-1, NB, 32 // GS, GS).mean(-1, keepdim=True)
    fine = torch.round(left).clamp(-(2 ** (u - 1)), 2 ** (u - 1) - 1)
    return ((coarse.reshape(-1, NB, 32 // GS, GS) + fine).reshape(-1, NB, 32) * grid).reshape(-1, D)


def _exact_attend(case, seed):
    B, T, Hq, Hkv, u = (case[k] for k in ("B", "T", "Hq", "Hkv", "u"))
    K, V = _keys_values(B, Hkv, case["ctx"] + T, seed)
    q, mask, lens = _attend_inputs(case, seed)
    G, H = Hq // Hkv, _hadamard64()
    sees = ((mask[:, :, None] >> torch.arange(T, device=DEV)) & 1).bool()
    out = torch.zeros((B, T, Hq, D), dtype=torch.float64, device=DEV)
    for b in range(B):
        n = int(lens[b])
        visible = torch.cat((torch.ones((T, n), dtype=torch.bool, device=DEV), sees[b]), 1)[:, None]
        for h in range(Hkv):
            k, v = _stored64(K[b, h, : n + T].double() @ H, u), _stored64(V[b, h, : n + T], u)
            s = (q[b, :, h * G:(h + 1) * G].double() @ H.T) @ k.T / math.sqrt(D)
            out[b, :, h * G:(h + 1) * G] = torch.softmax(s.masked_fill(~visible, -math.inf), -1) @ v
    return out


def _exact_write(case, seed):
    qkv, gain, _, start, pos, counts = _write_inputs(case, seed)
    B, T, Hq = case["B"], case["T"], case["Hq"]
    x = qkv.reshape(B, T, -1, D)[:, :, :Hq].double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * gain.double()
    at = (start[:, None] + torch.arange(T, device=DEV) if pos is None else pos).double()
    angle = at[..., None] / 500000.0 ** (torch.arange(0, D, 2, device=DEV).double() / D)
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    y = torch.view_as_real(torch.view_as_complex(y.reshape(B, T, Hq, D // 2, 2)) * turn).reshape(B, T, Hq, D)
    if counts is not None:
        y[torch.arange(T, device=DEV) >= counts[:, None]] = 0.0
    return [y] + [None] * 6


def exact(case, seed):
    """Verification and the move of rows give whole numbers only."""
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    return _exact_write(case, seed) if case["kind"] == "write" else None
