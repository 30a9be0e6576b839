"""The tree attention where a thread block walks many tiles of keys, and the verification where a warp walks many pieces of the
vocabulary: against plain forms in 64 bits on the GPU."""

import numpy as np
import pytest
import torch

from conftest import F32_REL_FRO_TOL
from oracle import tree_oracle as tro
from test_gpu_tree import _bf, _bound, _cache, _check_verify, _i32, _random_parents, _verify_case

pytestmark = pytest.mark.gpu

D = 128
RAGGED = [5900, 130, 260, 2000, 5, 383, 6000, 1400, 77, 3100]


def _gen(rng):
    return torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))


def _fields(plane, width, count):
    """Bytes [..., n] of a dense little-endian run of two's-complement fields -> float64 [..., count]."""
    bits = (plane[..., None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
    bits = bits.reshape(*plane.shape[:-1], -1)[..., :count * width].reshape(*plane.shape[:-1], count, width)
    weight = torch.tensor([2.0 ** k for k in range(width - 1)] + [-2.0 ** (width - 1)], dtype=torch.float64, device="cuda")
    return (bits.double() * weight).sum(-1)


def _values(planes, u):
    """Planes of gs = 2 with 32-blocks [Hkv, 4, L, ...] -> values [Hkv, L, 128] in 64 bits."""
    e, upper, shared = planes
    q = _fields(upper, 8 - u, 32) * 2.0 ** u + _fields(shared, u, 16).repeat_interleave(2, -1)
    x = q * torch.exp2(e.double())[..., None]
    return x.permute(0, 2, 1, 3).reshape(e.shape[0], e.shape[2], D)


def _hadamard():
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    while len(h) < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h / D ** 0.5


def _plain(q, c, lens, seen):
    """tro.tree_attention, one (sequence, kv head) at a time as matrices."""
    B, T, Hq, _ = q.shape
    G, H = Hq // c.Hkv, _hadamard()
    words = torch.from_numpy(np.stack([tro.mask_words(s) for s in seen])).cuda()
    sees = ((words[..., None] >> torch.arange(T, device="cuda")) & 1).bool()
    qd = torch.from_numpy(q).cuda().double()
    if c.rotate:
        qd = qd @ H
    out, mag, all_v = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(3))
    big = torch.zeros(q.shape[:3], dtype=torch.float64, device="cuda")
    for b in range(B):
        n = int(lens[b]) + T
        K, V = (_values([p[b, :, :, :n] for p in pl], c.u) for pl in (c.k, c.v))
        ok = torch.cat((torch.ones((T, n - T), dtype=torch.bool, device="cuda"), sees[b]), 1).repeat_interleave(G, 0)
        none = ~ok.any(1)
        for h in range(c.Hkv):
            x = qd[b, :, h * G:(h + 1) * G].reshape(T * G, D)
            s = (x @ K[h].T / D ** 0.5).masked_fill(~ok, -np.inf)
            p = torch.softmax(s.masked_fill(none[:, None], 0.0), -1).masked_fill(none[:, None], 0.0)
            a = (x.abs() @ K[h].abs().T / D ** 0.5).masked_fill(~ok, 0.0).amax(1)
            put = lambda t, y: t[b, :, h * G:(h + 1) * G].copy_(y.reshape(T, G, *y.shape[1:]))
            put(out, p @ V[h]), put(mag, p @ V[h].abs()), put(all_v, ok.double() @ V[h].abs()), put(big, a)
    return [t.cpu().numpy() for t in (out, mag, big, all_v)]


def _tiles(lens, T, Hkv, G):
    """Tiles of 128 keys of all items: row groups of 16, 32 or 64 rows."""
    R = T * G
    rows = 16 if R <= 16 else 32 if R <= 32 else 64
    return sum(-(-(int(n) + T) // 128) for n in lens) * Hkv * -(-R // rows)


def _case(rng, B, T, Hq, Hkv, u, lens, edit=None, aim=0.0, scale=1.0, least=4.0):
    """Fills a cache (keys along one direction per head, `aim` times how far into the context a key is) -> cache, queries, mask, lens,
    seen.  `least`: tiles per SM that the case has at least."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _tiles(lens, T, Hkv, Hq // Hkv) >= least * sms
    Lk = int(max(lens)) + T
    c = _cache(B, Hkv, D, (Lk + 15) // 16 * 16, u, 2, fill=0x7F)
    g = _gen(rng)
    w = torch.randn((1, Hkv, 1, D), generator=g, device="cuda")
    K, V = (torch.randn((B, Hkv, Lk, D), generator=g, device="cuda") for _ in range(2))
    K += aim * w * (torch.arange(Lk, device="cuda") / Lk)[:, None]
    q = torch.randn((B, T, Hkv, Hq // Hkv, D), generator=g, device="cuda") * scale
    if aim:
        q += w.reshape(Hkv, 1, D)
    if edit is not None:
        edit(K, V)
    for b in range(B):
        n = int(lens[b]) + T
        for X, pl, rot in ((K, c.k, True), (V, c.v, False)):
            part = [p[b:b + 1].contiguous() for p in pl]
            torch.ops.msaq.kv_write_into(X[b:b + 1, :, :n].to(torch.bfloat16).contiguous(), *part, Hkv, n, D, 4, 0, c.Lcap, u, 2, rot)
            for p, s in zip(pl, part):
                p[b:b + 1] = s
    seen = [tro.tree_mask(_random_parents(rng, T)) for _ in range(B)]
    mask = torch.from_numpy(np.stack([tro.mask_words(s) for s in seen])).cuda()
    q = q.reshape(B, T, Hq, D).to(torch.bfloat16).float().cpu().numpy()
    return c, q, mask, np.asarray(lens), seen


def _check(case, p_step=2.0 ** -11):
    c, q, mask, lens, seen = case
    Lk = int(max(lens)) + q.shape[1]
    got = c.attend_tree(_bf(q), mask, Lk, _i32(lens))
    again = c.attend_tree(_bf(q), mask, Lk, _i32(lens))
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    got = got.float().cpu().numpy()
    assert np.isfinite(got).all()
    ref, mag, big, all_v = _plain(q, c, lens, seen)
    err, lim = np.abs(got - ref), _bound(ref, mag, big, all_v, p_step)
    assert (err <= lim).all(), "worst %.3f of the bound" % (err / lim).max()
    return got, ref


# T and query heads to a kv head: 16, 32, 64 rows, and three groups of 64 of which the last is not full
ROWS = [(8, 2), (16, 2), (16, 4), (47, 3)]


@pytest.mark.parametrize("u", [4, 3, 2])
@pytest.mark.parametrize("T,G", ROWS)
def test_runs_of_many_tiles(rng, T, G, u):
    """Items longer and shorter than a run: ring slots, barriers and buffers are used again and again, queries of several items staged
    in one run, items finished in it or cut."""
    _check(_case(rng, 10, T, 8 * G, 8, u, RAGGED))


@pytest.mark.parametrize("aim", [1.5, 6.0, -3.0])
@pytest.mark.parametrize("T,G", ROWS)
def test_maximum_moves_within_a_run(rng, T, G, aim):
    """Scores that rise along the context (by 25 to 100 powers of two), or fall: references move while accumulators hold earlier tiles."""
    _check(_case(rng, 10, T, 8 * G, 8, 4, RAGGED, aim=aim, scale=0.3))


@pytest.mark.parametrize("u", [4, 2])
@pytest.mark.parametrize("T,G", ROWS)
def test_narrow_and_wide_values_in_a_run(rng, T, G, u):
    """Tiles whose values leave the range of fp16 between tiles whose values do not."""
    def edit(K, V):
        V[:, ::2, 300:310] *= 2.0 ** 12
        V[:, 1::2, 777] *= 2.0 ** 14
        V[:, :, 900:1100] *= 2.0 ** -26
        V[:, :, 2048:2050] *= 2.0 ** -40
        K[:, :, 512:640] *= 3

    _check(_case(rng, 10, T, 8 * G, 8, u, RAGGED, edit=edit), 2.0 ** -8)


@pytest.mark.parametrize("T,G", ROWS)
def test_batch_of_more_than_32_sequences(rng, T, G):
    """75 sequences of short, very short and no context; items of one tile beside items of several."""
    lens = rng.integers(0, 300, 75)
    lens[[3, 31, 32, 64, 70]] = [0, 128 - T, 129 - T, 0, 900]
    _check(_case(rng, 75, T, 4 * G, 4, 4, lens, least=2.0))


def test_few_long_sequences_cut_into_runs(rng):
    """Every item cut into many runs, some of which begin in the middle of one item and end in the middle of the next."""
    _check(_case(rng, 2, 8, 16, 8, 4, [9999, 6001]))


def _fp32(c, q, mask, Lk, lens):
    """The result before its rounding to bf16 (float32 output of the C ABI)."""
    from ms_kernel_b200 import _lib
    L, (B, T, Hq, _) = _lib.lib(), q.shape
    qd, ld = _bf(q), _i32(lens)
    out, of = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda"), torch.empty(q.shape, device="cuda")
    n = L.msaq_kv_tree_workspace(B, T, Hq, c.Hkv, Lk, D)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    _lib.check(L.msaq_kv_tree_attention(qd.data_ptr(), *[t.data_ptr() for t in (*c.k, *c.v)], out.data_ptr(), of.data_ptr(), ld.data_ptr(),
                                        mask.data_ptr(), T, B, T, Hq, c.Hkv, Lk, D, 4, c.u, c.gs, c.Lcap, 1, ws.data_ptr(), n,
                                        torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(of.to(torch.bfloat16), out)
    return of.double().cpu().numpy()


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("u", [4, 3, 2])
@pytest.mark.parametrize("T,G", ROWS)
def test_result_before_its_rounding(rng, T, G, u, far):
    """As near to 64 bits as the framework's other kernels before their rounding to bf16 (F32_REL_FRO_TOL), values far apart or not.
    Elementwise: a probability is held to 2^-20 of itself (2^-15 beside far values), a query element to 2^-21, sums to 2^-18, the
    smallest numbers of fp16 are 2^-31 of the largest probability."""
    def edit(K, V):
        V[:, ::2, ::300] *= 2.0 ** 12
        V[:, 1::2, 70::500] *= 2.0 ** -26

    c, q, mask, lens, seen = _case(rng, 10, T, 8 * G, 8, u, RAGGED, edit=edit if far else None)
    got = _fp32(c, q, mask, int(max(lens)) + T, lens)
    ref, mag, big, all_v = _plain(q, c, lens, seen)
    err, p = np.abs(got - ref), 2.0 ** -15 if far else 2.0 ** -20
    lim = mag * (2 * p + 2 * 2.0 ** -21 * big[..., None] + 2.0 ** -18 * (1 + big[..., None])) + 2.0 ** -31 * all_v
    assert np.linalg.norm(err) <= F32_REL_FRO_TOL * np.linalg.norm(ref)
    assert (err <= lim).all(), "worst %.3f of the bound" % (err / lim).max()


def _nodes_only(rng, u, gs, Lcap, T, ctx, K, V, seen, Hq=4):
    """One sequence, one kv head, given keys and values [ctx + T, 128] -> (result, reference, mag, big, all_v), fp32 and 64 bits."""
    c = _cache(1, 1, D, Lcap, u, gs, rotate=False)
    for X, pl in ((K, c.k), (V, c.v)):
        torch.ops.msaq.kv_write_into(X[None, None].to(torch.bfloat16).contiguous(), *pl, 1, ctx + T, D, 4, 0, Lcap, u, gs, False)
    q = np.zeros((1, T, Hq, D), np.float32)
    q[..., 0] = 1                                              # a key's first channel, over sqrt(128), is its score
    mask = torch.from_numpy(tro.mask_words(seen)).cuda()
    got = c.attend_tree(_bf(q), mask, ctx + T, _i32([ctx])).double().cpu().numpy()
    ref, mag, big, all_v = tro.tree_attention(q, [t.cpu().numpy() for t in c.k], [t.cpu().numpy() for t in c.v], u, gs, [ctx], [seen], False)
    return got, ref, mag, big, all_v


# the tuned kernel; another group size, another capacity: the generic one
KERNELS = [(4, 2, 0), (3, 2, 0), (2, 2, 0), (4, 8, 0), (4, 2, 1)]


@pytest.mark.parametrize("u,gs,odd", KERNELS)
@pytest.mark.parametrize("bits", [100, 110, 118, 120, 124, 126])
@pytest.mark.parametrize("ctx", [1, 4096])
def test_large_values_average_to_finite_numbers(rng, u, gs, odd, bits, ctx):
    """One key of 2^bits, or 4096 of them, and among the nodes one with a weight of 2^-30 and one of 2^-60 in front of them."""
    T, g = 4, _gen(rng)
    K, V = torch.zeros((ctx + T, D), device="cuda"), torch.ones((ctx + T, D), device="cuda")
    V[:ctx] *= 2.0 ** bits * (1 + 0.9 * torch.rand((ctx, D), generator=g, device="cuda"))
    V[ctx:] = torch.randn((T, D), generator=g, device="cuda").clamp(-3.9, 3.9)          # (times 2^126 still a number)
    V[ctx + 1] *= 2.0 ** bits
    K[ctx + 1, 0], K[ctx + 2, 0] = -235.0, -470.0              # e^(-235 / sqrt(128)) = 2^-30
    seen = [{0}, {0, 1}, {0, 2}, {3}]
    got, ref, mag, big, all_v = _nodes_only(rng, u, gs, (ctx + T + 15) // 16 * 16 + odd, T, ctx, K, V, seen)
    assert np.isfinite(got).all()
    err, lim = np.abs(got - ref), _bound(ref, mag, big, all_v, 2.0 ** -15)
    assert (err <= lim).all(), "worst %.3f of the bound" % (err / lim).max()


@pytest.mark.parametrize("u,gs,odd", KERNELS)
@pytest.mark.parametrize("bits", [110, 120, 126])
def test_small_values_beside_large_ones(rng, u, gs, odd, bits):
    """Nodes that attend only small values keep their digits beside nodes that attend large ones: a large value with a weight of 2^-30
    is a large number, the others are as if it were not there."""
    T, ctx, g = 6, 0, _gen(rng)
    K, V = torch.zeros((T, D), device="cuda"), torch.randn((T, D), generator=g, device="cuda")
    V[1] *= 2.0 ** -60
    V[3] = 2.0 ** bits * (1 + 0.9 * torch.rand(D, generator=g, device="cuda"))
    K[3, 0] = -235.0
    seen = [{0}, {1}, {0, 2}, {2, 3}, {4}, {1, 5}]
    got, ref, mag, big, all_v = _nodes_only(rng, u, gs, 16 + odd, T, ctx, K, V, seen)
    err, lim = np.abs(got - ref), _bound(ref, mag, big, all_v, 2.0 ** -15)
    assert (err <= lim).all(), "worst %.3f of the bound" % (err / lim).max()


@pytest.mark.parametrize("T,G", ROWS)
def test_large_values_in_a_run(rng, T, G):
    """Large values come up in the middle of some items, in front of and behind tiles of ordinary ones, while references move."""
    def edit(K, V):
        V[::2, ::3, 1500:1503] *= 2.0 ** 117
        V[1::2, 1::3, 64] *= 2.0 ** 121
        V[0, 2, 5000] *= 2.0 ** 95
        V[:, :, 200:210] *= 2.0 ** 13

    _check(_case(rng, 10, T, 8 * G, 8, 4, RAGGED, edit=edit, aim=2.0, scale=0.5), 2.0 ** -15)


@pytest.mark.parametrize("u", [4, 3, 2])
def test_values_without_a_finite_number(rng, u):
    """An infinity: NaN in the rows that attend it, the others as without it.  The largest finite values are numbers."""
    T, ctx = 5, 3
    for value in (2.0 ** 127, np.inf, -np.inf):
        K, V = torch.zeros((ctx + T, D), device="cuda"), torch.randn((ctx + T, D), generator=_gen(rng), device="cuda")
        V[ctx + 2, 77] = value
        seen = [{0}, {1}, {0, 2}, {2}, {0, 4}]
        c = _cache(1, 1, D, 16, u, 2, rotate=False)
        for X, pl in ((K, c.k), (V, c.v)):
            torch.ops.msaq.kv_write_into(X[None, None].to(torch.bfloat16).contiguous(), *pl, 1, ctx + T, D, 4, 0, 16, u, 2, False)
        q = _bf(rng.standard_normal((1, T, 4, D)))
        mask = torch.from_numpy(tro.mask_words(seen)).cuda()
        got = c.attend_tree(q, mask, ctx + T, _i32([ctx])).float().cpu().numpy()
        assert np.isfinite(got[0, [0, 1, 4]]).all()
        if np.isinf(value):
            assert np.isnan(got[0, 2:4]).all()
        else:
            assert np.isfinite(got).all()
        planes = [[t.cpu().numpy() for t in pl] for pl in (c.k, c.v)]
        planes[1][0][0, 0, :, ctx + 2] = 0                     # not attended by the others: any finite value will do
        ref, mag, big, all_v = tro.tree_attention(q.float().cpu().numpy(), *planes, u, 2, [ctx], [seen], False)
        ok = (np.abs(got - ref) <= _bound(ref, mag, big, all_v, 2.0 ** -15))[0, [0, 1, 4]]
        assert ok.all()


@pytest.mark.parametrize("bits", [-98, -95, -90])
def test_values_next_to_the_smallest_that_the_format_holds(rng, bits):
    """The quantiser's smallest block (2^-100 and below) counts as zeros; what is larger counts."""
    T, ctx = 2, 130
    K, V = torch.zeros((ctx + T, D), device="cuda"), 2.0 ** bits * (1 + 0.9 * torch.rand((ctx + T, D), generator=_gen(rng), device="cuda"))
    got, ref, mag, big, all_v = _nodes_only(rng, 4, 2, 144, T, ctx, K, V, [{0}, {0, 1}])
    lim = _bound(ref, mag, big, all_v, 2.0 ** -15) - 1e-30
    assert (np.abs(got - ref) <= lim).all()


@pytest.mark.parametrize("u,gs,odd", KERNELS)
@pytest.mark.parametrize("T,ctx", [(6, 45), (6, 126), (64, 100), (33, 0)])
def test_slots_that_nobody_attends_do_not_matter(rng, T, ctx, u, gs, odd):
    """Whatever bytes the slots hold that no mask bit names, inside the tree and behind it: the same bits come out."""
    B, Hq, Hkv, Lcap = 2, 8, 2, (ctx + T + 20) // 16 * 16 + odd
    c = _cache(B, Hkv, D, Lcap, u, gs)
    c.fill(*(_bf(rng.standard_normal((B, Hkv, ctx + T, D))) for _ in range(2)))
    parents = [[-1] + [0 if i % 3 else -1 for i in range(1, T)], [-1] * T]
    seen = [tro.tree_mask(p) for p in parents]
    seen[1][T - 1] = {0, T - 1}
    mask = torch.from_numpy(np.stack([tro.mask_words(s) for s in seen])).cuda()
    q, lens, outs = _bf(rng.standard_normal((B, T, Hq, D))), _i32([ctx, ctx - ctx // 3]), []
    for pattern in (None, 0x00, 0x7F, 0x80, 0x5A, 0xFF):
        if pattern is not None:
            for b in range(B):
                n = int(lens[b])
                free = sorted(set(range(T)) - set().union(*seen[b]))
                at = torch.tensor([n + j for j in free] + list(range(n + T, Lcap)), device="cuda")
                for t in (*c.k, *c.v):
                    t[b, :, :, at] = pattern - 256 if t.dtype == torch.int8 and pattern > 127 else pattern
        outs.append(c.attend_tree(q, mask, ctx + T, lens))
        assert torch.isfinite(outs[-1]).all() and torch.equal(outs[0], outs[-1]), pattern


@pytest.mark.parametrize("T,G", ROWS)
def test_rows_without_numbers_stay_alone_in_a_run(rng, T, G):
    """Queries with a NaN or an infinity: NaN in their rows, to the bit the same in all others."""
    c, q, mask, lens, _ = _case(rng, 10, T, 8 * G, 8, 4, RAGGED)
    Lk, ld = int(max(lens)) + T, _i32(lens)
    want = c.attend_tree(_bf(q), mask, Lk, ld)
    bad = torch.zeros(q.shape[:3], dtype=torch.bool)
    for b, i, h, d, x in ((0, 0, 0, 5, np.nan), (0, T - 1, 3, 0, np.inf), (4, 3, 8 * G - 1, 127, -np.inf), (6, 5, 1, 64, np.nan), (9, 2, 9, 1, np.inf)):
        q[b, i, h, d] = x
        bad[b, i, h] = True
    got = c.attend_tree(_bf(q), mask, Lk, ld)
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("stage", [0, 1, 4, 7])
@pytest.mark.parametrize("T,G,u", [(8, 2, 4), (16, 2, 3), (16, 4, 4), (47, 3, 2)])
def test_give_up_in_the_middle_of_a_run(rng, T, G, u, stage):
    """The first thread block's product of tile `stage` is never signalled: the items that its run touches are NaN, all others are as
    ever, the status word says so, and the next call is right."""
    import cabi
    c, q, mask, lens, _ = _case(rng, 10, T, 8 * G, 8, u, RAGGED, least=8.0)
    qd, ld, Lk = _bf(q), _i32(lens), int(max(lens)) + T
    want = c.attend_tree(qd, mask, Lk, ld)
    run = _tiles(lens, T, 8, G) // torch.cuda.get_device_properties(0).multi_processor_count
    assert run > stage
    torch.ops.msaq.wait_status(True)
    with cabi.options({3: 4096, 4: stage}):
        got = c.attend_tree(qd, mask, Lk, ld)
        torch.cuda.synchronize()
    assert torch.ops.msaq.wait_status(True) == 4
    R, tile = T * G, 0
    rows = 16 if R <= 16 else 32 if R <= 32 else 64
    for b in range(len(lens)):
        for hk in range(8):
            x, y = (t[b, :, hk * G:(hk + 1) * G].reshape(R, D) for t in (got, want))
            for r0 in range(0, R, rows):
                if tile < run:
                    assert torch.isnan(x[r0:r0 + rows]).all(), (b, hk, r0)
                else:
                    assert torch.equal(x[r0:r0 + rows], y[r0:r0 + rows]), (b, hk, r0)
                tile += -(-(int(lens[b]) + T) // 128)
    assert torch.equal(c.attend_tree(qd, mask, Lk, ld), want)
    assert torch.ops.msaq.wait_status(True) == 0


# ------------------------------------------------------------------------------------------------ verify_tree
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V,dtype", [(65536, torch.float32), (65537, torch.float32), (70001, torch.bfloat16), (128256, torch.float32),
                                     (200003, torch.bfloat16)])
def test_verify_large_vocabularies(rng, V, dtype, drawn):
    """More than 512 entries to a warp."""
    p, d, tokens, parents, u = _verify_case(rng, 3, 6, V, drawn, near=2.0)
    parents[0, 1:] = 0                                         # a chain of rejections
    _check_verify(p, d, tokens, parents, u, dtype)
