"""CPU checks of the operators of a step with several drafted tokens: refusals before anything touches a device, the tree helper, and
the oracle's own properties."""

import numpy as np
import pytest
import torch

from oracle import tree_oracle as tro


def test_write_qkv_refuses():
    from ms_kernel_b200 import _lib
    L, one = _lib.lib(), 16

    def call(**kw):
        a = dict(qkv=one, ld=1536, q=one, k=[one] * 3, v=[one] * 3, B=2, T=3, H=8, Hkv=2, D=128, NB=4, start=0, sp=None, pos=None, counts=None,
                 qg=one, kg=one, f32=0, eps=1e-6, cos=one, sin=one, rows=64, Lcap=64, u=4, gs=2, rot=1)
        a.update(kw)
        return L.msaq_kv_write_qkv(a["qkv"], a["ld"], a["q"], *a["k"], *a["v"], a["B"], a["T"], a["H"], a["Hkv"], a["D"], a["NB"], a["start"],
                                   a["sp"], a["pos"], a["counts"], a["qg"], a["kg"], a["f32"], a["eps"], a["cos"], a["sin"], a["rows"],
                                   a["Lcap"], a["u"], a["gs"], a["rot"], None)

    for bad in (dict(qkv=None), dict(q=None), dict(k=[one, None, one]), dict(B=0), dict(T=0), dict(Hkv=-1), dict(NB=3), dict(ld=1535),
                dict(start=62), dict(start=-1), dict(cos=None), dict(sin=None), dict(rows=1), dict(rows=2), dict(sp=one, rows=63),
                dict(eps=-1.0), dict(eps=float("nan")), dict(k=[one, one + 1, one]), dict(f32=1, qg=one + 2), dict(B=1 << 20, T=1 << 20, Lcap=1 << 21)):
        assert call(**bad) == -1, bad
    for bad in (dict(D=96, NB=3, ld=4096), dict(u=5), dict(gs=3)):
        assert call(**bad) == -2, bad
    if not torch.cuda.is_available():
        assert call() == -5 and call(cos=None, sin=None, rows=0) == -5 and call(T=1, rows=1) == -5 and call(pos=one, rows=2) == -5


def test_tree_attention_refuses():
    from ms_kernel_b200 import _lib
    L, one = _lib.lib(), 16

    def call(**kw):
        a = dict(q=one, k=[one] * 3, v=[one] * 3, out=one, mask=one, stride=0, B=2, T=8, H=8, Hkv=2, Lk=64, D=128, NB=4, u=4, gs=2, Lcap=64, ws=one,
                 wsb=1 << 40)
        a.update(kw)
        return L.msaq_kv_tree_attention(a["q"], *a["k"], *a["v"], a["out"], None, None, a["mask"], a["stride"], a["B"], a["T"], a["H"], a["Hkv"],
                                        a["Lk"], a["D"], a["NB"], a["u"], a["gs"], a["Lcap"], 1, a["ws"], a["wsb"], None)

    for bad in (dict(q=None), dict(mask=None), dict(out=None), dict(v=[one, one, None]), dict(T=0), dict(T=65), dict(B=0), dict(H=9), dict(NB=2),
                dict(Lk=7), dict(Lcap=63), dict(stride=7), dict(mask=20), dict(k=[one, 18, one]), dict(B=65536), dict(H=1 << 20, Hkv=1 << 20)):
        assert call(**bad) == -1, bad
    for bad in (dict(D=48), dict(u=1), dict(gs=64)):
        assert call(**bad) == -2, bad
    assert L.msaq_kv_tree_workspace(0, 8, 8, 2, 64, 128) == 0 and L.msaq_kv_tree_workspace(1, 65, 8, 2, 128, 128) == 0
    assert L.msaq_kv_tree_workspace(1, 8, 8, 2, 64, 128) > 65536
    if not torch.cuda.is_available():
        assert call() == -5


def test_verify_and_keep_refuse():
    from ms_kernel_b200 import _lib
    L, one = _lib.lib(), 16

    def verify(**kw):
        a = dict(p=one, psb=800, pst=100, q=None, qsb=0, qst=0, f32=1, tok=one, par=one, parsb=0, u=one, path=one, count=one, token=one, B=2, T=8, V=100)
        a.update(kw)
        return L.msaq_verify_tree(a["p"], a["psb"], a["pst"], a["q"], a["qsb"], a["qst"], a["f32"], a["tok"], a["par"], a["parsb"], a["u"],
                                  a["path"], a["count"], a["token"], a["B"], a["T"], a["V"], None)

    for bad in (dict(p=None), dict(tok=None), dict(u=None), dict(token=None), dict(B=0), dict(T=0), dict(T=65), dict(V=0), dict(V=(1 << 30) + 1),
                dict(psb=-1), dict(q=one, qst=-1), dict(p=18), dict(q=17, f32=0)):
        assert verify(**bad) == -1, bad

    def keep(**kw):
        a = dict(k=[one] * 3, v=[one] * 3, path=one, count=one, start=0, sp=None, B=2, T=8, Hkv=2, NB=4, Lcap=64, u=4, gs=2)
        a.update(kw)
        return L.msaq_kv_keep(*a["k"], *a["v"], a["path"], a["count"], a["start"], a["sp"], a["B"], a["T"], a["Hkv"], a["NB"], a["Lcap"], a["u"],
                              a["gs"], None)

    for bad in (dict(path=None), dict(count=None), dict(k=[None, one, one]), dict(T=65), dict(T=0), dict(B=0), dict(start=57), dict(start=-1),
                dict(v=[one, 18, one]), dict(B=1 << 30)):
        assert keep(**bad) == -1, bad
    assert keep(u=7) == -2
    if not torch.cuda.is_available():
        assert verify() == -5 and keep() == -5


def test_operators_refuse_cpu_tensors():
    from ms_kernel_b200 import ops
    p = torch.rand(1, 2, 8)
    i = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.verify_tree(p, i, i, torch.rand(1, 2))
    cache = ops.KVCache(1, 2, 128, 32, 4, 2, "cpu")
    with pytest.raises(RuntimeError):
        cache.write_qkv(torch.zeros(1, 2, 8 * 128, dtype=torch.bfloat16), 4, 0)
    with pytest.raises(RuntimeError):
        cache.attend_tree(torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16), torch.ones(2, dtype=torch.int64), 8)
    with pytest.raises(RuntimeError):
        cache.keep(0, i, torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        cache.keep(0, torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        cache.attend_tree(torch.zeros(2, 2, 4, 128, dtype=torch.bfloat16), torch.ones(2, dtype=torch.int64), 8)


def test_write_qkv_refuses_another_batch_than_the_cache():
    from ms_kernel_b200 import ops
    cache = ops.KVCache(3, 2, 128, 32, 4, 2, "cpu")
    for B in (2, 4):
        with pytest.raises(ValueError):
            cache.write_qkv(torch.zeros(B, 1, 8 * 128, dtype=torch.bfloat16), 4, 0)


def test_tree_attention_refuses_more_keys_than_its_indexes_hold():
    from ms_kernel_b200 import _lib
    L, one, most = _lib.lib(), 16, 1 << 30

    def call(Lk):
        return L.msaq_kv_tree_attention(one, *[one] * 3, *[one] * 3, one, None, None, one, 0, 1, 8, 1, 1, Lk, 32, 1, 4, 2, (1 << 31) - 1, 1, one,
                                        1 << 40, None)

    assert L.msaq_kv_tree_workspace(1, 8, 1, 1, most, 32) > 65536 and L.msaq_kv_tree_workspace(1, 8, 1, 1, most + 1, 32) == 0
    assert call(most + 1) == -1
    if not torch.cuda.is_available():
        assert call(most) == -5


@pytest.mark.parametrize("T", [1, 2, 7, 64])
def test_tree_mask_against_sets(rng, T):
    from ms_kernel_b200 import ops
    rows = []
    for _ in range(3):
        par = [-1] + [int(rng.integers(-1, i)) for i in range(1, T)]
        rows.append(par)
    mask, depth = ops.tree_mask(rows, "cpu")
    assert mask.dtype == torch.int64 and depth.dtype == torch.int32 and tuple(mask.shape) == (3, T)
    for b, par in enumerate(rows):
        seen = tro.tree_mask(par)
        assert np.array_equal(mask[b].numpy(), tro.mask_words(seen))
        assert [max(len(s) - 1, 0) for s in seen] == depth[b].tolist()
    m1, d1 = ops.tree_mask(np.array(rows[0]), "cpu")
    assert torch.equal(m1, mask[0]) and torch.equal(d1, depth[0])


def test_tree_mask_refuses():
    from ms_kernel_b200 import ops
    for bad in ([0, 0], [-1, 1], [-1, 0, 3], [-1, -2], [], np.zeros((1, 2, 2), int), [-1] + list(range(64))):
        with pytest.raises(ValueError):
            ops.tree_mask(bad, "cpu")


@pytest.mark.parametrize("drawn", [False, True])
def test_oracle_verification_keeps_the_targets_distribution(drawn):
    """The first token behind the root has the target's distribution, whatever the drafts: frequencies of 40000 steps over a vocabulary
    of five, each within five standard deviations (below 0.0125)."""
    rng = np.random.default_rng(5)
    V, n = 5, 40000
    p = np.array([0.4, 0.25, 0.2, 0.1, 0.05])
    q = np.array([0.1, 0.3, 0.15, 0.2, 0.25])
    target, draft = np.tile(p, (4, 1)), np.tile(q, (4, 1))
    got = np.zeros(V)
    for _ in range(n):
        toks = rng.choice(V, 3, p=q) if drawn else np.array([1, 0, 4])
        tokens = np.concatenate([[0], toks])
        path, token = tro.verify_tree(target, tokens, [-1, 0, 0, 0], rng.random(4), draft if drawn else None)
        got[tokens[path[1]] if len(path) > 1 else token] += 1
    assert np.abs(got / n - p).max() < 0.0125


def test_tree_attention_refuses_a_workspace_that_is_not_aligned():
    """Partial results are read sixteen bytes at a time."""
    from ms_kernel_b200 import _lib
    L, one = _lib.lib(), 16

    def call(ws):
        return L.msaq_kv_tree_attention(one, *[one] * 3, *[one] * 3, one, None, None, one, 0, 1, 8, 8, 2, 64, 128, 4, 4, 2, 64, 1, ws, 1 << 40, None)

    for ws in (one + 1, one + 4, one + 8):
        assert call(ws) == -1
    if not torch.cuda.is_available():
        assert call(one) == -5 and call(None) == -5


def test_write_qkv_refuses_positions_of_another_shape():
    """[T, B] has as many elements as [B, T]: taken as it stands, it would give most tokens another token's position."""
    from ms_kernel_b200 import ops
    cache = ops.KVCache(2, 2, 128, 32, 4, 2, "cpu")
    qkv = torch.zeros(2, 3, 8 * 128, dtype=torch.bfloat16)
    for shape in ((3, 2), (1, 6), (2, 4)):
        with pytest.raises(ValueError):
            cache.write_qkv(qkv, 4, 0, pos=torch.zeros(shape, dtype=torch.int32))
    with pytest.raises(RuntimeError):                          # this one is only on the wrong device
        cache.write_qkv(qkv, 4, 0, pos=torch.zeros(2, 3, dtype=torch.int32))


def test_tree_mask_refuses_a_number():
    from ms_kernel_b200 import ops
    with pytest.raises(ValueError):
        ops.tree_mask(-1, "cpu")
