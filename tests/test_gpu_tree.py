"""GPU parity of the operators of a step with several drafted tokens against their plain forms in 64 bits."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import msaq_oracle as orc
from oracle import tree_oracle as tro

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _bf(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16).cuda()


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _planes(planes):
    return [t.cpu().numpy() for t in planes]


def _status(clear=True):
    return torch.ops.msaq.wait_status(clear)


def _random_parents(rng, T):
    return [-1] + [int(i - 1 if rng.random() < 0.5 else rng.integers(0, i)) for i in range(1, T)]


def _cache(B, Hkv, D, Lcap, u, gs, rotate=True, fill=None):
    from ms_kernel_b200 import ops
    c = ops.KVCache(B, Hkv, D, Lcap, u, gs, "cuda", rotate=rotate)
    if fill is not None:
        for t in (*c.k, *c.v):
            t.fill_(fill if t.dtype == torch.int8 else fill & 0xFF)
    return c


# ------------------------------------------------------------------------------------------------ write_qkv
def _check_write(rng, B, T, Hq, Hkv, D, u, gs, Lcap, rotate=True, gains="bf16", rope=True, start=None, pos=None, counts=None, slack=0):
    c = _cache(B, Hkv, D, Lcap, u, gs, rotate, fill=0x5A)
    width = (Hq + 2 * Hkv) * D
    qkv = orc.to_bf16(rng.standard_normal((B, T, width)).astype(np.float32) * rng.uniform(0.2, 3, (1, 1, width)).astype(np.float32))
    dev = torch.zeros((B * T, width + slack), dtype=torch.bfloat16, device="cuda")
    dev[:, :width] = _bf(qkv.reshape(B * T, width))
    x = torch.as_strided(dev, (B, T, width), (T * (width + slack), width + slack, 1))
    start = rng.integers(0, Lcap - T + 1, B) if start is None else start
    g = [None, None]
    if gains:
        g = [1 + 0.3 * rng.standard_normal(D).astype(np.float32) for _ in range(2)]
        g = [orc.to_bf16(a) for a in g] if gains == "bf16" else g
    gd = [None if a is None else (_bf(a) if gains == "bf16" else torch.from_numpy(a).cuda()) for a in g]
    tables = orc.rope_tables(np.arange(Lcap), D) if rope else None
    td = None if tables is None else tuple(torch.from_numpy(t).cuda() for t in tables)
    pk, pv = _planes(c.k), _planes(c.v)
    want = tro.write_qkv(qkv, pk, pv, Hq, Hkv, D, u, gs, start, tables, g[0], g[1], EPS, pos, counts, rotate)
    q = c.write_qkv(x, Hq, _i32(start), td, gd[0], gd[1], EPS, pos=None if pos is None else _i32(pos),
                    counts=None if counts is None else _i32(counts))
    assert tuple(q.shape) == (B, T, Hq, D) and q.dtype == torch.bfloat16
    assert np.array_equal(q.float().cpu().numpy(), want)
    for got, ref in zip((*c.k, *c.v), (*pk, *pv)):
        assert np.array_equal(got.cpu().numpy(), ref)


@pytest.mark.parametrize("u,gs", [(4, 2), (3, 2), (2, 2), (4, 8), (3, 4), (2, 32)])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_write_every_format_and_head_dim(rng, u, gs, D):
    _check_write(rng, 2, 5, 6, 2, D, u, gs, 23)


@pytest.mark.parametrize("B,T,Hq,Hkv", [(1, 1, 32, 8), (1, 1, 1, 1), (3, 1, 7, 7), (1, 61, 8, 1), (2, 33, 5, 1), (1, 130, 12, 4)])
def test_write_heads_and_lengths(rng, B, T, Hq, Hkv):
    _check_write(rng, B, T, Hq, Hkv, 128, 4, 2, T + 9)


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("gains", [None, "bf16", "fp32"])
@pytest.mark.parametrize("rope", [False, True])
def test_write_with_and_without_norm_rope_rotation(rng, rotate, gains, rope):
    _check_write(rng, 2, 4, 4, 2, 128, 4, 2, 16, rotate=rotate, gains=gains, rope=rope)
    _check_write(rng, 2, 4, 4, 2, 64, 3, 4, 16, rotate=rotate, gains=gains, rope=rope)


@pytest.mark.parametrize("u,gs", [(4, 2), (4, 4)])
def test_write_trees_padding_and_strides(rng, u, gs):
    B, T, Lcap = 3, 6, 40
    start = rng.integers(0, 20, B)
    pos = start[:, None] + np.array([[0, 1, 1, 2, 2, 3]])
    counts = np.array([6, 1, 0])
    for slack in (0, 8, 3):                                    # 3: rows that are not 16-byte aligned
        _check_write(rng, B, T, 4, 2, 128, u, gs, Lcap, start=start, pos=pos, counts=counts, slack=slack)


def test_write_skips_and_reports_what_is_outside(rng):
    _status()
    Lcap, T = 12, 4
    _check_write(rng, 3, T, 4, 2, 128, 4, 2, Lcap, start=np.array([-2, 3, 10]))
    assert _status() == 8
    _check_write(rng, 2, T, 4, 2, 128, 4, 8, Lcap, start=np.array([9, -1]))
    assert _status() == 8
    pos = np.array([[0, 1, -1, 3], [4, 12, 6, 7]])
    _check_write(rng, 2, T, 4, 2, 128, 4, 2, Lcap, start=np.array([0, 4]), pos=pos)
    assert _status() == 8
    _check_write(rng, 2, T, 4, 2, 128, 4, 2, Lcap, start=np.array([0, 4]))
    assert _status() == 0


def test_write_equals_the_append_of_one_token(rng):
    """Without a norm a token's bytes are those of append with RoPE."""
    B, Hq, Hkv, D, Lcap, at = 2, 8, 2, 128, 32, 17
    qkv = _bf(rng.standard_normal((B, 1, (Hq + 2 * Hkv) * D)))
    tables = tuple(torch.from_numpy(t).cuda() for t in orc.rope_tables(np.arange(Lcap), D))
    a, b = _cache(B, Hkv, D, Lcap, 4, 2), _cache(B, Hkv, D, Lcap, 4, 2)
    q = a.write_qkv(qkv, Hq, at, tables)
    heads = qkv.reshape(B, Hq + 2 * Hkv, D)
    b.append(heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:], at, tables)
    for x, y in zip((*a.k, *a.v), (*b.k, *b.v)):
        assert torch.equal(x, y)
    one = tuple(t[at:at + 1].contiguous() for t in tables)
    assert torch.equal(q[:, 0], torch.ops.msaq.rope(heads[:, :Hq].contiguous(), *one, None, 0))


def test_write_norm_of_extreme_rows(rng):
    """Zero rows, rows whose squares leave the range of fp32, one huge channel."""
    Hq, Hkv, D, Lcap = 4, 1, 128, 16
    c = _cache(1, Hkv, D, Lcap, 4, 2)
    x = rng.standard_normal((1, 1, Hq + 2 * Hkv, D)).astype(np.float32)
    x[0, 0, 0] = 0
    x[0, 0, 1] *= 1e30
    x[0, 0, 2] *= 1e-30
    x[0, 0, 3, 7] = 1e20
    x[0, 0, 4] *= 1e25
    x = orc.to_bf16(x)
    g = orc.to_bf16(1 + 0.3 * rng.standard_normal(D).astype(np.float32))
    pk, pv = _planes(c.k), _planes(c.v)
    want = tro.write_qkv(x.reshape(1, 1, -1), pk, pv, Hq, Hkv, D, 4, 2, [3], None, g, g, EPS, None, None, True)
    q = c.write_qkv(_bf(x.reshape(1, 1, -1)), Hq, 3, None, _bf(g), _bf(g), EPS)
    assert np.array_equal(q.float().cpu().numpy(), want)
    for got, ref in zip((*c.k, *c.v), (*pk, *pv)):
        assert np.array_equal(got.cpu().numpy(), ref)


@pytest.mark.parametrize("T,Hq,Hkv,D,u", [(2601, 10, 3, 128, 4), (4321, 10, 3, 128, 4), (7201, 10, 3, 128, 3), (7201, 9, 5, 64, 2), (1999, 40, 9, 256, 4),
                                            (1500, 10, 3, 128, 4), (800, 10, 3, 128, 2), (400, 10, 3, 128, 3)])
def test_write_prompt_equals_its_pieces(rng, T, Hq, Hkv, D, u):
    """A long prompt (several heads in a row per lane, the last run shorter) writes what its pieces of 97 tokens write one by one,
    to the bit, with two sequences, padding, positions that are not the slots and tables on a 4-byte boundary."""
    B, Lcap = 2, T + 40
    qkv = _bf(rng.standard_normal((B, T, (Hq + 2 * Hkv) * D), dtype=np.float32))
    gains = [_bf(1 + 0.3 * rng.standard_normal(D)) for _ in range(2)]
    tables = [torch.from_numpy(t).cuda() for t in orc.rope_tables(np.arange(Lcap), D)]
    moved = [torch.cat([t.new_zeros(1), t.flatten()])[1:].view_as(t) for t in tables]
    assert moved[0].data_ptr() % 16 == 4
    start, counts = np.array([3, 17]), np.array([T, T - 111])
    pos = (np.arange(T)[None] // 2 + start[:, None]).astype(np.int32)
    a, b = _cache(B, Hkv, D, Lcap, u, 2, fill=0x5A), _cache(B, Hkv, D, Lcap, u, 2, fill=0x5A)
    q = a.write_qkv(qkv, Hq, _i32(start), tables, *gains, EPS, pos=_i32(pos), counts=_i32(counts))
    for t in range(0, T, 97):
        n = min(97, T - t)
        part = b.write_qkv(qkv[:, t:t + n].contiguous(), Hq, _i32(start + t), moved, *gains, EPS, pos=_i32(pos[:, t:t + n]),
                           counts=_i32(np.clip(counts - t, 0, n)))
        assert torch.equal(part, q[:, t:t + n])
    for x, y in zip((*a.k, *a.v), (*b.k, *b.v)):
        assert torch.equal(x, y)
    assert _status() == 0


# ------------------------------------------------------------------------------------------------ attend_tree
def _bound(ref, mag, big, all_v, p_step):
    """Elementwise bound of the output's error, relative steps of half a unit: the result's rounding to bf16 (2^-8 of it); of a
    probability (p_step: 2^-11 in fp16, 2^-8 in bf16) and, twice -- numerator and denominator --, what a score is off by: a
    query element is held in fp16 at least (2^-11), which moves a score by 2^-11 sum |q_d k_d| / sqrt(D) at most; and 2^-18 for sums in 32 bits.
    fp16 ends: its smallest number is 2^-24, so a probability held times 2^7 relative to the largest one (or to one up to 2^8 smaller) is
    off by up to 2^-25 / 2^7 = 2^-32 of the largest, whatever its own size; the largest is at most the sum of all, so the average moves by
    2^-32 sum |v| at most."""
    return 2.0 ** -8 * np.abs(ref) + mag * (2 * p_step + 2 * 2.0 ** -11 * big[..., None] + 2.0 ** -18 * (1 + big[..., None])) + 2.0 ** -32 * all_v + 1e-30


def _attend_case(rng, B, T, Hq, Hkv, D, u, gs, lens, Lcap, rotate=True, seen=None, shared=False, scale=1.0, edit=None, p_step=2.0 ** -11):
    c = _cache(B, Hkv, D, Lcap, u, gs, rotate, fill=0x7F)      # slots that nothing names hold the largest exponent
    Lk = int(max(lens)) + T
    K = orc.to_bf16(rng.standard_normal((B, Hkv, Lk, D)).astype(np.float32) * scale)
    V = orc.to_bf16(rng.standard_normal((B, Hkv, Lk, D)).astype(np.float32))
    if edit is not None:
        edit(K, V)
    kd, vd = _bf(K), _bf(V)
    for b in range(B):                                         # only what a sequence has; the rest stays as it was
        n = int(lens[b]) + T
        for X, pl, rot in ((kd, c.k, rotate), (vd, c.v, False)):
            part = [p[b:b + 1].contiguous() for p in pl]
            torch.ops.msaq.kv_write_into(X[b:b + 1, :, :n].contiguous(), *part, Hkv, n, D, D // 32, 0, Lcap, u, gs, rot)
            for p, s in zip(pl, part):
                p[b:b + 1] = s
    if seen is None:
        seen = [tro.tree_mask(_random_parents(rng, T)) for _ in range(B)]
        if shared:
            seen = [seen[0]] * B
    words = np.stack([tro.mask_words(s) for s in seen])
    mask = torch.from_numpy(words[0] if shared else words).cuda()
    q = orc.to_bf16(rng.standard_normal((B, T, Hq, D)).astype(np.float32) * scale)
    got = c.attend_tree(_bf(q), mask, Lk, _i32(lens)).float().cpu().numpy()
    ref, mag, big, all_v = tro.tree_attention(q, _planes(c.k), _planes(c.v), u, gs, lens, seen, rotate)
    assert np.isfinite(got).all()
    err = np.abs(got - ref)
    lim = _bound(ref, mag, big, all_v, p_step)
    assert (err <= lim).all(), "worst %.3f of the bound" % (err / lim).max()
    return c, q, mask, Lk, got


FORMATS = [(4, 2), (3, 2), (2, 2), (4, 8), (3, 16), (2, 4)]


@pytest.mark.parametrize("u,gs", FORMATS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_attend_every_format_and_head_dim(rng, u, gs, D):
    _attend_case(rng, 2, 5, 6, 2, D, u, gs, np.array([37, 150]), 160)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (8, 2), (6, 2), (10, 2), (7, 1), (8, 1), (12, 1), (32, 8)])
@pytest.mark.parametrize("T", [1, 8, 13])
def test_attend_heads(rng, Hq, Hkv, T):
    _attend_case(rng, 1, T, Hq, Hkv, 128, 4, 2, np.array([131]), 160)


@pytest.mark.parametrize("u", [4, 3, 2])
@pytest.mark.parametrize("T", [1, 2, 3, 16, 17, 31, 33, 63, 64])
def test_attend_tree_sizes(rng, T, u):
    _attend_case(rng, 2, T, 4, 1, 128, u, 2, np.array([100, 61]), 208)


@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 17, 111, 112, 127, 128, 129, 255, 1000])
def test_attend_context_lengths(rng, ctx):
    _attend_case(rng, 1, 9, 4, 2, 128, 4, 2, np.array([ctx]), (ctx + 9 + 15) // 16 * 16)


@pytest.mark.parametrize("u", [4, 3])
def test_attend_long_ragged_batch(rng, u):
    _attend_case(rng, 4, 6, 8, 2, 128, u, 2, np.array([2500, 0, 1203, 2047]), 2512)


@pytest.mark.parametrize("rotate", [False, True])
def test_attend_capacity_and_shared_tree(rng, rotate):
    _attend_case(rng, 2, 7, 8, 2, 128, 4, 2, np.array([90, 33]), 101, rotate=rotate, shared=True)   # capacity no multiple of 16
    _attend_case(rng, 2, 7, 8, 2, 128, 4, 2, np.array([90, 33]), 112, rotate=rotate, shared=True)


@pytest.mark.parametrize("u,gs", [(4, 2), (4, 8)])
def test_attend_masks_that_leave_rows_empty(rng, u, gs):
    """No context and no node named: zeros; a row that names others but not itself; bits beyond the tree count for nothing."""
    T = 6
    seen = [[set(), {0}, {0, 2}, {5}, {1, 3}, {0, 63, 40}], [set(), set(), {2}, {0, 1, 2}, {4}, {1}]]
    _, _, _, _, got = _attend_case(rng, 2, T, 8, 2, 128, u, gs, np.array([0, 19]), 32, seen=seen)
    assert (got[0, 0] == 0).all()


@pytest.mark.parametrize("u,gs", [(4, 2), (3, 2), (4, 8)])
def test_attend_infinities_in_unseen_nodes(rng, u, gs):
    """A node whose key and value are infinite or NaN in the model reaches only the rows that attend it."""
    B, T, Hq, Hkv, D, lens, Lcap = 1, 6, 8, 2, 128, np.array([45]), 64
    bad = 3
    seen = [[{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 2, 4}, {0, 5}]]

    def edit(K, V):
        K[:, :, 45 + bad], V[:, :, 45 + bad] = np.inf, -np.inf
        V[:, :, 45 + bad, ::3] = np.nan

    c = _cache(B, Hkv, D, Lcap, u, gs, fill=0x7F)
    n = 45 + T
    K = rng.standard_normal((B, Hkv, n, D)).astype(np.float32)
    V = rng.standard_normal((B, Hkv, n, D)).astype(np.float32)
    edit(K, V)
    c.fill(_bf(K), _bf(V))
    q = orc.to_bf16(rng.standard_normal((B, T, Hq, D)).astype(np.float32))
    mask = torch.from_numpy(np.stack([tro.mask_words(s) for s in seen])).cuda()
    got = c.attend_tree(_bf(q), mask, n, _i32(lens)).float().cpu().numpy()
    rows = [i for i in range(T) if bad not in seen[0][i]]
    pk, pv = _planes(c.k), _planes(c.v)
    for pl in (*pk, *pv):
        pl[:, :, :, 45 + bad] = 0                              # not attended by these rows: any finite value will do
    keep = [[s if bad not in s else set() for s in seen[0]]]
    ref, mag, big, all_v = tro.tree_attention(q, pk, pv, u, gs, lens, keep, True)
    lim = _bound(ref, mag, big, all_v, 2.0 ** -8)
    assert np.isfinite(got[:, rows]).all()
    assert (np.abs(got - ref)[:, rows] <= lim[:, rows]).all()


@pytest.mark.parametrize("u", [4, 3, 2])
def test_attend_value_ranges_far_apart(rng, u):
    """Value rows of 2^-90 to 2^90 in one tile, seen by different nodes: no row loses its digits to another's range."""
    T = 5
    seen = [[{0}, {1}, {2}, {3}, {0, 3}]]
    scales = [2.0 ** -90, 2.0 ** -30, 1.0, 2.0 ** 90, 2.0 ** -60]

    def edit(K, V):
        for i in range(T):
            V[:, :, i] *= scales[i]

    _attend_case(rng, 1, T, 4, 1, 128, u, 2, np.array([0]), 16, seen=seen, edit=edit, p_step=2.0 ** -8)


def test_attend_key_ranges_far_apart(rng):
    """Keys of very different size, and query rows of very different size, in one call."""
    def edit(K, V):
        K[:, :, ::3] *= 2.0 ** -40
        K[:, :, 1::7] *= 16

    _attend_case(rng, 1, 8, 8, 2, 128, 4, 2, np.array([200]), 208, edit=edit)


def test_attend_dominant_key_far_in_front(rng):
    """One key far above all others early on: later tiles weigh next to nothing, and the other way round."""
    for at in (3, 600):
        def edit(K, V):
            K[:, :, at] *= 12
        _attend_case(rng, 1, 8, 4, 1, 128, 4, 2, np.array([900]), 912, edit=edit, scale=1.5)


def test_attend_nan_query_row_stays_alone(rng):
    c, q, mask, Lk, got = _attend_case(rng, 1, 8, 8, 2, 128, 4, 2, np.array([70]), 80)
    q2 = q.copy()
    q2[0, 3, 5, 17] = np.nan
    q2[0, 6, 0, 99] = np.inf
    again = c.attend_tree(_bf(q2), mask, Lk, _i32([70])).float().cpu().numpy()
    assert np.isnan(again[0, 3, 5]).all() and np.isnan(again[0, 6, 0]).all()
    same = np.ones(got.shape, bool)
    same[0, 3, 5] = same[0, 6, 0] = False
    assert np.array_equal(again[same], got[same])


def test_attend_one_node_is_ordinary_decoding(rng):
    """T = 1 attends what attend attends: both within the bound, and lens clipped to the cache's keys."""
    c, q, mask, Lk, got = _attend_case(rng, 2, 1, 8, 2, 128, 4, 2, np.array([99, 40]), 112)
    plain = c.attend(_bf(q)[:, 0], Lk, _i32([100, 41])).float().cpu().numpy()
    assert orc.rel_fro(got[:, 0], plain) < 2.0 ** -7
    far = c.attend_tree(_bf(q), mask, Lk, _i32([5000, -3]))     # clipped to Lk - T and to 0
    near = c.attend_tree(_bf(q), mask, Lk, _i32([99, 0]))
    assert torch.equal(far, near)
    full, named = c.attend_tree(_bf(q), mask, Lk), c.attend_tree(_bf(q), mask, Lk, _i32([99, 99]))
    assert torch.equal(full[0], named[0])                       # (the second sequence's slots from 41 on stand for no numbers)


def test_attend_fp32_output_is_what_is_rounded(rng):
    from ms_kernel_b200 import _lib
    c, q, mask, Lk, got = _attend_case(rng, 1, 8, 8, 2, 128, 4, 2, np.array([300]), 320)
    L = _lib.lib()
    qd, out, of = _bf(q), torch.empty(q.shape, dtype=torch.bfloat16, device="cuda"), torch.empty(q.shape, device="cuda")
    n = L.msaq_kv_tree_workspace(1, 8, 8, 2, Lk, 128)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    args = [qd.data_ptr(), *[t.data_ptr() for t in (*c.k, *c.v)], out.data_ptr(), of.data_ptr(), None, mask.data_ptr(), 8, 1, 8, 8, 2, Lk, 128, 4,
            4, 2, c.Lcap, 1, ws.data_ptr()]
    assert L.msaq_kv_tree_attention(*args, n - 1, None) == -3
    _lib.check(L.msaq_kv_tree_attention(*args, n, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(of.to(torch.bfloat16), out) and np.array_equal(out.float().cpu().numpy(), got)


# ------------------------------------------------------------------------------------------------ verify_tree
def _softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _verify_case(rng, B, T, V, drawn, near=1.0, shared=False):
    z = rng.standard_normal((B, T, V)) * 2
    p = _softmax(z)
    d = _softmax(z + near * rng.standard_normal((B, T, V)))
    parents = np.array([_random_parents(rng, T) for _ in range(B)], np.int32)
    if shared:
        parents[:] = parents[0]
    tokens = np.zeros((B, T), np.int32)
    for b in range(B):
        for j in range(1, T):
            row = d[b, parents[b, j]].astype(np.float64)
            tokens[b, j] = rng.choice(V, p=row / row.sum()) if drawn else int(np.argsort(-row, kind="stable")[(parents[b, :j] == parents[b, j]).sum() % V])
    return p, (d if drawn else None), tokens, parents, rng.random((B, T)).astype(np.float32)


def _check_verify(p, d, tokens, parents, u, dtype=torch.float32, shared=False):
    from ms_kernel_b200 import ops
    pt = torch.from_numpy(p).cuda().to(dtype)
    dt = None if d is None else torch.from_numpy(d).cuda().to(dtype)
    par = torch.from_numpy(parents[0] if shared else parents).cuda()
    path, count, token = ops.verify_tree(pt, torch.from_numpy(tokens).cuda(), par, torch.from_numpy(u).cuda(), dt)
    pn = pt.float().cpu().numpy()
    dn = None if d is None else dt.float().cpu().numpy()
    lengths = []
    for b in range(len(p)):
        want, tok = tro.verify_tree(pn[b], tokens[b], parents[b], u[b], None if dn is None else dn[b])
        assert path[b].tolist() == want + [-1] * (p.shape[1] - len(want)), b
        assert int(count[b]) == len(want) and int(token[b]) == tok, b
        lengths.append(len(want))
    return lengths


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (2, 2, 2), (5, 9, 3), (3, 16, 127), (4, 33, 128), (2, 64, 1001), (3, 8, 4096), (2, 12, 32003)])
def test_verify_against_the_plain_form(rng, B, T, V, drawn):
    _check_verify(*_verify_case(rng, B, T, V, drawn))


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("near", [0.0, 5.0])
def test_verify_drafts_equal_and_far(rng, drawn, near):
    """Drafts drawn from the target itself are all accepted on a chain; far ones reject again and again."""
    p, d, tokens, parents, u = _verify_case(rng, 4, 20, 500, drawn, near)
    if drawn and near == 0.0:
        parents[:] = np.arange(20) - 1
        d = p.copy()
        for b in range(4):
            for j in range(1, 20):
                tokens[b, j] = rng.choice(500, p=p[b, j - 1].astype(np.float64) / p[b, j - 1].sum(dtype=np.float64))
        assert _check_verify(p, d, tokens, parents, u) == [20] * 4
    else:
        _check_verify(p, d, tokens, parents, u)


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_bf16_probabilities_and_shared_tree(rng, drawn):
    p, d, tokens, parents, u = _verify_case(rng, 3, 12, 777, drawn, shared=True)
    _check_verify(p, d, tokens, parents, u, torch.bfloat16, shared=True)
    _check_verify(p, d, tokens, parents, u, torch.float32, shared=True)


def test_verify_siblings_with_one_token_and_nodes_that_are_not_there(rng):
    p, d, tokens, parents, u = _verify_case(rng, 6, 16, 50, True, near=3.0)
    parents[:, 1:] = 0
    tokens[:, 4] = tokens[:, 3]
    parents[1, 5:] = -1
    parents[2, 6] = 9                                          # not in front of it
    tokens[3, 2:6] = [-1, 50, 1 << 30, -(1 << 31)]             # outside the vocabulary
    parents[4, 3] = 1 << 30
    for drafts in (d, None):
        _check_verify(p, drafts, tokens, parents, u)


def test_verify_empty_infinite_and_negative_probabilities(rng):
    p, d, tokens, parents, u = _verify_case(rng, 6, 8, 300, True)
    p[0, :] = 0                                                # nothing anywhere: no token
    p[1, 0] = d[1, 0]                                          # nothing left of p after a rejection
    p[1, 0, tokens[1, 1]] = 0
    p[2, :, ::5] = np.nan
    p[3, :, 1::4] = -1
    p[4, :, 2::9] = np.inf
    d[5, :, ::3] = np.nan
    u[1] = 0.999
    for drafts in (d, None):
        _check_verify(p, drafts, tokens, parents, u)


def test_verify_greedy_targets_and_edges_of_the_draw(rng):
    """One-hot targets follow the drafts exactly; random numbers 0 and just below 1; tokens without probability are never drawn."""
    B, T, V = 4, 6, 1000
    p = np.zeros((B, T, V), np.float32)
    best = rng.integers(0, V, (B, T))
    for b in range(B):
        for i in range(T):
            p[b, i, best[b, i]] = 1
    parents = np.tile(np.arange(T, dtype=np.int32) - 1, (B, 1))
    tokens = np.zeros((B, T), np.int32)
    tokens[:, 1:] = best[:, :-1]
    tokens[1, 3] = (tokens[1, 3] + 1) % V                       # wrong from its third node on
    u = np.zeros((B, T), np.float32)
    u[2:] = np.nextafter(np.float32(1), np.float32(0))
    assert _check_verify(p, None, tokens, parents, u) == [6, 3, 6, 6]
    q = _softmax(rng.standard_normal((B, T, V)))
    q[:, :, 100:] = 0
    _check_verify(q, None, tokens, parents, u)


def test_verify_strided_rows(rng):
    from ms_kernel_b200 import ops
    p, d, tokens, parents, u = _verify_case(rng, 3, 7, 130, True)
    want = ops.verify_tree(*(torch.from_numpy(x).cuda() for x in (p, tokens, parents, u, d)))
    for pad in (1, 4):
        wide = torch.full((3, 9, 130 + pad), 7.0, device="cuda")
        wide[:, 1:8, pad:] = torch.from_numpy(p).cuda()
        dr = torch.full((7, 3, 130 + pad), 7.0, device="cuda")
        dr[:, :, :130] = torch.from_numpy(d).cuda().transpose(0, 1)
        got = ops.verify_tree(wide[:, 1:8, pad:], *(torch.from_numpy(x).cuda() for x in (tokens, parents, u)), dr.transpose(0, 1)[..., :130])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ keep
@pytest.mark.parametrize("u,gs,D", [(4, 2, 128), (3, 2, 128), (2, 2, 64), (4, 8, 32), (3, 32, 256), (2, 16, 128)])
@pytest.mark.parametrize("T", [1, 7, 33, 64])
def test_keep_moves_the_accepted_rows(rng, u, gs, D, T):
    B, Hkv, Lcap = 4, 3, T + 21
    c = _cache(B, Hkv, D, Lcap, u, gs)
    for t in (*c.k, *c.v):
        t.copy_(torch.randint(0, 127, t.shape, device="cuda").to(t.dtype))
    start = rng.integers(0, Lcap - T + 1, B)
    path = np.full((B, T), -1, np.int32)
    count = np.zeros(B, np.int32)
    for b in range(B):
        way = sorted(rng.choice(T, int(rng.integers(1, T + 1)), replace=False)) if b else []
        path[b, :len(way)], count[b] = way, len(way)
    if T > 2:
        path[3, :3], count[3] = [2, 0, 2], 3                   # any order, a node twice
    want = [tro.keep(_planes(pl), start, path, count) for pl in (c.k, c.v)]
    c.keep(_i32(start), _i32(path), _i32(count))
    for pl, ref in zip((c.k, c.v), want):
        for got, r in zip(pl, ref):
            assert np.array_equal(got.cpu().numpy(), r)
    assert _status() == 0


def test_keep_skips_and_reports_what_is_outside(rng):
    _status()
    B, T, Lcap = 3, 4, 16
    c = _cache(B, 2, 128, Lcap, 4, 2)
    c.fill(_bf(rng.standard_normal((B, 2, Lcap, 128))), _bf(rng.standard_normal((B, 2, Lcap, 128))))
    before = [t.clone() for t in (*c.k, *c.v)]
    c.keep(_i32([-1, 14, 0]), _i32([[1, 2, 3, -1], [3, 3, -1, -1], [4, -2, 1 << 30, 0]]), _i32([3, 2, 3]))
    assert _status() == 8
    for a, b in zip(before, (*c.k, *c.v)):
        assert torch.equal(a, b)
    c.keep(0, _i32([[0, 1, 2, 3]] * B), _i32([9, -5, 0]))       # counts beyond the path are clipped
    assert _status() == 0
    for a, b in zip(before, (*c.k, *c.v)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ together
class _ToyModel:
    """Embedding -> QKV of a token, one attention layer, probabilities of the next token."""

    def __init__(self, rng, V, Hq, Hkv, D, Lcap):
        self.V, self.Hq, self.Hkv, self.D = V, Hq, Hkv, D
        self.table = _bf(rng.standard_normal((V, (Hq + 2 * Hkv) * D)))
        self.head = torch.from_numpy(rng.standard_normal((Hq * D, V)).astype(np.float32) * 0.3).cuda()
        self.rope = tuple(torch.from_numpy(t).cuda() for t in orc.rope_tables(np.arange(Lcap), D))
        self.qg, self.kg = (_bf(1 + 0.2 * rng.standard_normal(D)) for _ in range(2))

    def nodes(self, cache, tokens, mask, lens, depth, Lk):
        """tokens int32 [B,T] -> probabilities [B,T,V]; the nodes' keys and values are in the cache then."""
        qkv = self.table[tokens.long()]
        q = cache.write_qkv(qkv, self.Hq, lens, self.rope, self.qg, self.kg, EPS, pos=(lens[:, None] + depth).to(torch.int32))
        a = cache.attend_tree(q, mask, Lk, lens)
        return torch.softmax(a.reshape(*tokens.shape, -1).float() @ self.head, -1), a


@pytest.mark.parametrize("u,gs", [(4, 2), (3, 2), (4, 8)])
def test_speculative_steps_leave_the_cache_of_plain_decoding(rng, u, gs):
    """Write, attend, verify, keep over several steps; then the accepted tokens one at a time through another cache: the
    same bytes in every slot in front of the root, and the last node's attention alike."""
    from ms_kernel_b200 import ops
    B, T, V, Hq, Hkv, D, Lcap, steps = 3, 7, 40, 8, 2, 128, 128, 6
    m = _ToyModel(rng, V, Hq, Hkv, D, Lcap)
    par = [-1, 0, 0, 1, 1, 2, 3]
    mask, depth = ops.tree_mask(par)
    parents = _i32(par)
    cache = _cache(B, Hkv, D, Lcap, u, gs)
    prompt = rng.integers(0, V, (B, 5))
    counts = np.array([5, 3, 4])                               # a padded batch of prompts
    first = m.table[torch.from_numpy(prompt).cuda()]
    cache.write_qkv(first, Hq, 0, m.rope, m.qg, m.kg, EPS, counts=_i32(counts))
    lens = _i32(counts)
    history = [list(prompt[b, :counts[b]]) for b in range(B)]
    root = _i32(rng.integers(0, V, B))
    for _ in range(steps):
        tokens = _i32(rng.integers(0, V, (B, T)))
        tokens[:, 0] = root
        probs, _ = m.nodes(cache, tokens, mask, lens, depth, Lcap)
        probs = probs ** 0.2                                   # flatter, so that random drafts are accepted now and then
        probs = probs / probs.sum(-1, keepdim=True)
        path, count, token = ops.verify_tree(probs, tokens, parents, torch.from_numpy(rng.random((B, T)).astype(np.float32) * 0.05).cuda())
        cache.keep(lens, path, count)
        for b in range(B):
            history[b] += [int(tokens[b, i]) for i in path[b].tolist() if i >= 0]
        lens = lens + count
        root = token
    assert max(len(h) for h in history) > 5 + steps            # something was accepted
    other = _cache(B, Hkv, D, Lcap, u, gs)
    one_mask, one_depth = ops.tree_mask([-1])
    n = max(len(h) for h in history)
    for t in range(n):
        tok = _i32([[h[min(t, len(h) - 1)]] for h in history])
        at = _i32([min(t, len(h) - 1) for h in history])       # a shorter sequence writes its last token again
        _, a = m.nodes(other, tok, one_mask, at, one_depth.reshape(1, 1), Lcap)
    for b, h in enumerate(history):
        assert int(lens[b]) == len(h)
        for x, y in zip((*cache.k, *cache.v), (*other.k, *other.v)):
            assert torch.equal(x[b, :, :, :len(h)], y[b, :, :, :len(h)])


def test_steps_captured_and_replayed(rng):
    """The four calls in one CUDA graph: replays follow the lengths, tokens and probabilities in device memory."""
    from ms_kernel_b200 import ops
    B, T, V, Hq, Hkv, D, Lcap = 2, 5, 64, 8, 2, 128, 96
    m = _ToyModel(rng, V, Hq, Hkv, D, Lcap)
    par = [-1, 0, 0, 1, 2]
    mask, depth = ops.tree_mask(par)
    parents = _i32(par)
    runs = []
    for captured in (False, True):
        g = np.random.default_rng(3)
        cache = _cache(B, Hkv, D, Lcap, 4, 2)
        lens, root = _i32([11, 4]), _i32(g.integers(0, V, B))
        cache.write_qkv(m.table[torch.from_numpy(g.integers(0, V, (B, 11))).cuda()], Hq, 0, m.rope, m.qg, m.kg, EPS)
        tokens, u = torch.zeros((B, T), dtype=torch.int32, device="cuda"), torch.zeros((B, T), device="cuda")

        def step():
            probs, a = m.nodes(cache, tokens, mask, lens, depth, Lcap)
            path, count, token = ops.verify_tree(probs, tokens, parents, u)
            cache.keep(lens, path, count)
            lens.add_(count)
            tokens[:, 0] = token
            return path, a

        if captured:
            keep_state = [t.clone() for t in (lens, tokens, u, *cache.k, *cache.v)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = step()
            for t, s in zip((lens, tokens, u, *cache.k, *cache.v), keep_state):
                t.copy_(s)
        tokens[:, 0] = root
        log = []
        for _ in range(5):
            tokens[:, 1:] = torch.from_numpy(g.integers(0, V, (B, T - 1))).to(torch.int32).cuda()
            u.copy_(torch.from_numpy(g.random((B, T)).astype(np.float32) * 0.02))
            if captured:
                graph.replay()
                path, a = outs
            else:
                path, a = step()
            log += [path.clone(), a.clone(), lens.clone()]
        runs.append(log + [t.clone() for t in (*cache.k, *cache.v)])
    for x, y in zip(*runs):
        assert torch.equal(x, y)


def test_calls_on_two_streams_do_not_meet(rng):
    """The same calls on two streams at once, each with its own cache: the results of one after the other."""
    from ms_kernel_b200 import ops
    jobs = []
    for i in range(2):
        c, q, mask, Lk, got = _attend_case(rng, 1, 16, 8, 2, 128, 4, 2, np.array([1500 + i]), 1520)
        jobs.append((c, _bf(q), mask, Lk, got))
    p, d, tokens, parents, u = (torch.from_numpy(x).cuda() for x in _verify_case(rng, 4, 16, 5000, True))
    want = ops.verify_tree(p, tokens, parents, u, d)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(20):
        for s, (c, q, mask, Lk, _) in zip(streams, jobs):
            with torch.cuda.stream(s):
                outs.append((c.attend_tree(q, mask, Lk, None), ops.verify_tree(p, tokens, parents, u, d)))
    torch.cuda.synchronize()
    for i, (a, v) in enumerate(outs):
        assert np.array_equal(a.float().cpu().numpy(), jobs[i % 2][4])
        assert all(torch.equal(x, y) for x, y in zip(v, want))


def test_attend_gives_up_and_recovers(rng):
    """A product whose completion is never signalled: the waits run out, the rows are NaN, the status word says so, and the next call is
    right."""
    import cabi
    c, q, mask, Lk, got = _attend_case(rng, 1, 8, 8, 1, 128, 4, 2, np.array([1000]), 1008)
    _status()
    with cabi.options({3: 4096, 4: 0}):
        bad = c.attend_tree(_bf(q), mask, Lk)
        torch.cuda.synchronize()
    assert _status() == 4
    assert torch.isnan(bad).all()
    assert np.array_equal(c.attend_tree(_bf(q), mask, Lk).float().cpu().numpy(), got)
    assert _status() == 0
